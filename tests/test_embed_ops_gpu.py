"""Token embedding with its gradient by sorted ids (ops/csrc/embed_kernels.hip via
models/train_ops.py) against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _ref(ids, table, add, scale, dx):
    """x, dtable and sum |terms| of dtable, in 64 bits."""
    V, H = table.shape
    i, d = ids.reshape(-1).long(), dx.reshape(-1, H).double() * scale
    x = table.double()[i]
    g, mag = (torch.zeros(V, H, dtype=torch.float64, device=table.device) for _ in range(2))
    g.index_add_(0, i, d)
    mag.index_add_(0, i, d.abs())
    if add is not None:
        a = add.reshape(-1).long()
        at = a[a >= 0]
        x[a >= 0] += table.double()[at]
        g.index_add_(0, at, d[a >= 0])
        mag.index_add_(0, at, d[a >= 0].abs())
    return (x * scale).reshape(*ids.shape, H), g, mag


def _check(ids, table, add, scale, seed=0):
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(seed)
    t = table.dtype
    dx = torch.randn(*ids.shape, table.shape[1], generator=g, device=dev).to(t)
    leaf = table.detach().clone().requires_grad_()
    x = train_ops.embed_lookup(ids, leaf, add, scale=scale)
    (dt,) = torch.autograd.grad(x, leaf, dx)
    # the kernel takes the scale in fp32: so does the reference
    rx, rg, mag = _ref(ids, table, add, float(torch.tensor(scale, dtype=torch.float32)), dx)
    assert x.dtype == t and x.shape == (*ids.shape, table.shape[1]) and dt.dtype == t and dt.shape == table.shape
    # x: one sum, one product in fp32 and one rounding to the type; fp16 below its normal
    # range has a step of 2^-24 (half: 2^-25)
    tiny = 2.0 ** -25 if t == torch.float16 else 0.0
    two = 2 * 2.0 ** -24
    ax = (table.double().abs()[ids.long()] + (0 if add is None else
          table.double().abs()[add.long().clamp(min=0)] * (add >= 0).unsqueeze(-1))) * abs(scale)
    assert ((x.double() - rx).abs() <= rx.abs() * HALF_STEP[t] * 1.01 + ax * two + tiny).all()
    # dtable: n terms summed in fp32 (at most n roundings of at most sum |terms| each, in
    # practice far fewer in a tree of depth 64 + 4 + n / 64), the scale, and one to the type
    n = 2 * ids.numel() + 2
    depth = min(n, 64 + 64 + n // 64 + 8)
    assert ((dt.double() - rg).abs() <= rg.abs() * HALF_STEP[t] * 1.01 + mag * depth * 2.0 ** -24 + tiny).all()
    return x, dt


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,V,H", [(1, 1, 1), (45, 8192, 256), (128, 300, 65), (129, 5, 8), (257, 77, 96), (4001, 1000, 576),
                                   (8192, 40, 100), (8193, 8576, 64), (20011, 300000, 24),
                                   (300001, 500, 8)])
def test_embed_matches_definition(dtype, n, V, H):
    """Both sides of every rule: one launch / sort by ranges / radix passes, one to three 8-bit
    passes, 16-byte rows and odd ones, with and without a second row."""
    g = torch.Generator(device=dev).manual_seed(n)
    table = torch.randn(V, H, generator=g, device=dev).to(dtype)
    ids = torch.randint(0, V, (n,), generator=g, device=dev)
    add = torch.randint(-2, V, (n,), generator=g, device=dev)
    _check(ids, table, None, 1.0)
    _check(ids.int(), table, add.int(), 3.0 ** 0.5, seed=1)


@pytest.mark.parametrize("n", [200, 3000, 16000, 40000])
def test_embed_same_id_everywhere(n):
    """One id for every position (and a lone other at each end): the long-run path."""
    table = torch.randn(50, 72, device=dev)
    ids = torch.full((n,), 7, device=dev)
    ids[0], ids[-1] = 49, 0
    _check(ids, table, None, 1.0)
    _check(ids, table, torch.full((n,), 7, device=dev), 0.5)


def test_embed_repeats_bit_for_bit_and_takes_views():
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(3)
    table = torch.randn(600, 576, generator=g, device=dev)
    ids = torch.randint(0, 600, (61, 128), generator=g, device=dev).t()  # not contiguous
    x, dt = _check(ids, table, None, 1.0)
    for _ in range(3):
        x2, dt2 = _check(ids, table, None, 1.0)
        assert torch.equal(x, x2) and torch.equal(dt, dt2)
    # rows of a wider matrix (not contiguous), a table that starts off a 16-byte border
    wide = torch.randn(600, 70, generator=g, device=dev)
    _check(ids, wide[:, 3:68], None, 1.0)
    flat = torch.randn(600 * 64 + 1, generator=g, device=dev)
    _check(ids, flat[1:].view(600, 64), None, 1.0)
    # a gradient that autograd expands from one number
    leaf = table.clone().requires_grad_()
    train_ops.embed_lookup(ids, leaf).sum().backward()
    want = torch.zeros(600, device=dev).index_add_(0, ids.reshape(-1), torch.ones(ids.numel(), device=dev))
    assert torch.equal(leaf.grad, want[:, None].expand(-1, 576))


def test_embed_edges():
    """No ids at all; ids of no row: NaN, and nothing of them in the gradient."""
    from smsgate_amd.models import train_ops

    table = torch.randn(10, 8, device=dev, requires_grad=True)
    x = train_ops.embed_lookup(torch.empty(0, 3, dtype=torch.long, device=dev), table)
    assert x.shape == (0, 3, 8)
    assert not torch.autograd.grad(x.sum(), table)[0].any()
    for n in (5, 300, 17000):
        ids = torch.arange(n, device=dev) % 10
        bad = torch.arange(n, device=dev) % 5 == 4
        ids[bad] = torch.where(torch.arange(int(bad.sum()), device=dev) % 2 == 0, 10, -1)
        add = torch.full_like(ids, -7)
        x = train_ops.embed_lookup(ids, table, add)
        assert x[bad].isnan().all() and torch.equal(x[~bad], table[ids[~bad]])
        (dt,) = torch.autograd.grad(x, table, torch.ones_like(x))
        want = torch.zeros(10, device=dev).index_add_(0, ids[~bad], torch.ones(int((~bad).sum()), device=dev))
        assert torch.equal(dt, want[:, None].expand(-1, 8))
        far = torch.full_like(ids, 10)
        assert train_ops.embed_lookup(torch.zeros_like(ids), table, far).isnan().all()


def test_embed_streams_and_graph():
    """On a stream of its own, and captured: replays between eager calls on other ids."""
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(5)
    for n in (100, 5000, 20000):
        table = torch.randn(9000, 64, generator=g, device=dev)
        dx = torch.randn(n, 64, generator=g, device=dev)
        ids = torch.randint(0, 9000, (n,), generator=g, device=dev)

        def step(leaf):
            x = train_ops.embed_lookup(ids, leaf)
            return x, torch.autograd.grad(x, leaf, dx)[0]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            leaf = table.clone().requires_grad_()
            step(leaf)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gx, gd = step(leaf)
        for k in range(4):
            ids.copy_(torch.randint(0, 9000, (n,), generator=g, device=dev))
            want_x, want_d = step(table.clone().requires_grad_())
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(gx, want_x) and torch.equal(gd, want_d), (n, k)
