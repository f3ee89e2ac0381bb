"""The training operators (models/train_ops.py) where indexes pass 32 bits, where calls share
or repeat what they should not, and where ignored rows hold anything."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"


def test_embed_offsets_past_32_bits():
    """2.3e9 elements of x and dx: rows from both ends, and a gradient of ones (counts, exact)."""
    from smsgate_amd.models import train_ops

    n, V, H = 4_000_003, 777, 576
    ids = (torch.arange(n, device=dev) * 31) % V
    table = torch.randn(V, H, device=dev, requires_grad=True)
    x = train_ops.embed_lookup(ids, table)
    for s in (slice(0, 1000), slice(n // 2, n // 2 + 1000), slice(n - 1000, n)):
        assert torch.equal(x[s], table[ids[s]])
    (dt,) = torch.autograd.grad(x, table, torch.ones(1, device=dev).expand(n, H))
    want = torch.bincount(ids, minlength=V).float()
    assert torch.equal(dt, want[:, None].expand(-1, H))


def test_attention_offsets_past_32_bits():
    """4.4e9 elements of q (heads far apart in memory): a short sequence in a long, wide batch
    gives what it gives alone."""
    from smsgate_amd.models import train_ops

    nh, nkv, T, D, n = 520, 130, 131_072, 64, 100
    g = torch.Generator(device=dev).manual_seed(1)
    lengths = torch.tensor([n], dtype=torch.int32, device=dev)
    small = [torch.randn(1, h, n, D, generator=g, device=dev).bfloat16() for h in (nh, nkv, nkv)]
    dsmall = torch.randn(1, n, nh * D, generator=g, device=dev).bfloat16()
    far = []
    for t in small:
        big = torch.zeros(1, t.shape[1], T, D, dtype=torch.bfloat16, device=dev)
        big[:, :, :n] = t
        far.append(big.requires_grad_())
    dout = torch.zeros(1, T, nh * D, dtype=torch.bfloat16, device=dev)
    dout[:, :n] = dsmall
    near = [t.requires_grad_() for t in small]
    a = train_ops.tiled_attention(*near)
    want = torch.autograd.grad(a, near, dsmall)
    b = train_ops.tiled_attention(*far, lengths=lengths)
    assert torch.equal(b[:, :n], a) and not b[:, n:].any()
    got = torch.autograd.grad(b, far, dout)
    for x, y in zip(got, want):
        # one block of keys per key head here, one per query head in the short call: the
        # heads' sums may round apart by a step of the type
        assert float((x[:, :, :n].double() - y.double()).norm()) <= 2.0 ** -8 * float(y.double().norm())
        assert not x[:, :, n:].any()


def test_loss_offsets_past_32_bits():
    """2.3e9 elements of the table and its gradient, in eight pieces of the vocabulary."""
    from smsgate_amd.models import train_ops

    V, H, N = 4_000_003, 576, 5
    g = torch.Generator(device=dev).manual_seed(2)
    table = torch.empty(V, H, dtype=torch.bfloat16, device=dev)
    table.normal_(0.0, 0.05, generator=g)
    h = torch.randn(N, H, generator=g, device=dev).bfloat16()
    labels = torch.tensor([0, V - 1, V // 2, 7, V - 1], device=dev)
    h.requires_grad_(), table.requires_grad_()
    loss = train_ops.lm_loss(h, table, labels, reduction="sum")
    dh, dt = torch.autograd.grad(loss, (h, table))
    with torch.no_grad():
        step = 250_000
        x = h.double()
        z = torch.cat([x @ table[i:i + step].double().t() for i in range(0, V, step)], 1)
        lse = torch.logsumexp(z, 1)
        # 16 roundings of values up to 20 in each of 5 rows
        assert abs(float(loss) - float((lse - z.gather(1, labels[:, None])[:, 0]).sum())) <= 5 * 16 * 20 * 2.0 ** -24
        d = torch.exp(z - lse[:, None])
        d[torch.arange(N, device=dev), labels] -= 1.0
        want = sum(d[:, i:i + step] @ table[i:i + step].double() for i in range(0, V, step))
        assert float((dh.double() - want).norm()) <= 2 * 2.0 ** -8 * float(want.norm())
        for i in (0, V // 2 - 10, V - step):
            w = d[:, i:i + step].t() @ x
            assert float((dt[i:i + step].double() - w).norm()) <= 2 * 2.0 ** -8 * float(w.norm())


def test_ignored_rows_may_hold_anything():
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(3)
    h = torch.randn(300, 64, generator=g, device=dev).bfloat16()
    table = torch.randn(500, 64, generator=g, device=dev).bfloat16().requires_grad_()
    labels = torch.randint(0, 500, (300,), generator=g, device=dev)
    labels[::3] = -100
    dirty = h.clone()
    dirty[0::6], dirty[3::6] = math.nan, math.inf
    res = []
    for x in (h, dirty):
        x = x.requires_grad_()
        loss = train_ops.lm_loss(x, table, labels)
        res.append((loss.detach(), *torch.autograd.grad(loss, (x, table))))
    for a, b in zip(*res):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_one_key_has_no_gradient(dtype, causal):
    """A row that sees one key: P = 1, so dq and dk are 0, not what rounding leaves of dP - D."""
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(6)
    for T, lens in ((1, None), (70, [1, 1, 0]), (200, [1, 1, 1])):
        q, k, v = (torch.randn(3, h, T, 64, generator=g, device=dev).to(dtype).requires_grad_() for h in (6, 2, 2))
        lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
        out = train_ops.tiled_attention(q, k, v, causal=causal, lengths=lengths)
        dq, dk, dv = torch.autograd.grad(out, (q, k, v), torch.randn(out.shape, generator=g, device=dev).to(dtype))
        assert not dq.any() and not dk.any() and dv.any()
        n = 1 if lens is None else lens[0]
        assert torch.equal(out[0, :n].reshape(n, 6, 64), v[0, :, :n].transpose(0, 1).repeat_interleave(3, 1))
    q, k, v = (torch.randn(1, h, 100, 64, generator=g, device=dev).to(dtype).requires_grad_() for h in (6, 2, 2))
    out = train_ops.tiled_attention(q, k, v)
    (dq,) = torch.autograd.grad(out, q, torch.ones_like(out))
    assert not dq[:, :, 0].any() and dq[:, :, 1].any()


def test_sure_rows_lose_nothing():
    """The label's logit far above all others (or alone): the loss and the gradients are 0."""
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(8)
    for V, N in ((1, 5), (600, 200), (9000, 2100)):
        table = torch.randn(V, 64, generator=g, device=dev)
        table = (table / table.norm(dim=1, keepdim=True)).bfloat16()
        labels = torch.randint(0, V, (N,), generator=g, device=dev)
        h = (table[labels].float() * 900).bfloat16().requires_grad_()  # ahead by 900 (1 - cos)
        table.requires_grad_()
        each = train_ops.lm_loss(h, table, labels, reduction="none")
        far = (h.double() @ table.double().t()).topk(min(2, V), 1).values
        sure = torch.ones(N, dtype=torch.bool, device=dev) if V == 1 else far[:, 0] - far[:, 1] > 110.0
        assert sure.float().mean() > 0.9
        assert not each[sure].any()
        dh, dt = torch.autograd.grad(each, (h, table), sure.float())
        assert not dh.any() and not dt.any()


def _calls():
    """(name, leaves, a call of them) of each operator, small enough to be launched together."""
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(4)

    def normal(*s):
        return torch.randn(*s, generator=g, device=dev)

    ids = torch.randint(0, 900, (3000,), generator=g, device=dev)
    labels = torch.randint(-1, 900, (700,), generator=g, device=dev)
    lengths = torch.tensor([150, 80], dtype=torch.int32, device=dev)
    return [
        ("embed", [normal(900, 64).requires_grad_()], lambda t: train_ops.embed_lookup(ids, t)),
        ("attention", [normal(2, h, 150, 64).bfloat16().requires_grad_() for h in (6, 2, 2)],
         lambda q, k, v: train_ops.tiled_attention(q, k, v, lengths=lengths)),
        ("loss", [normal(700, 64).bfloat16().requires_grad_(), normal(900, 64).bfloat16().requires_grad_()],
         lambda h, t: train_ops.lm_loss(h, t, labels, reduction="none", ignore_index=-1)),
    ]


def test_backward_twice_gives_the_same():
    for name, leaves, call in _calls():
        out = call(*leaves)
        g = torch.ones_like(out)
        a = torch.autograd.grad(out, leaves, g, retain_graph=True)
        b = torch.autograd.grad(out, leaves, g)
        for x, y in zip(a, b):
            assert torch.equal(x, y), name


def test_no_second_derivatives():
    """Refused, not wrong."""
    for name, leaves, call in _calls():
        out = call(*leaves)
        grads = torch.autograd.grad(out, leaves, torch.ones_like(out).requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError):
            grads[0].float().sum().backward()


def test_calls_on_streams_at_once_do_not_meet():
    """The same calls on four streams, launched without waiting, against one at a time."""
    calls = _calls()
    want = []
    for name, leaves, call in calls:
        out = call(*leaves)
        want.append((out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                for name, leaves, call in calls:
                    out = call(*leaves)
                    got.append((name, (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))))
    torch.cuda.synchronize()
    for i, (name, res) in enumerate(got):
        for x, y in zip(res, want[i % len(calls)]):
            assert torch.equal(x, y), (name, i)
    del got


def test_two_graphs_of_one_pool():
    """Two captured graphs that share a memory pool, replayed in turn between eager calls."""
    calls = _calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs, pool = [], [], None
    with torch.cuda.stream(side):
        for name, leaves, call in calls:
            out = call(*leaves)
            torch.autograd.grad(out, leaves, torch.ones_like(out))
            del out  # no eager graph of the leaves lives while one is captured
    torch.cuda.current_stream().wait_stream(side)
    for name, leaves, call in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = call(*leaves)
            res = (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))
            del out
        graphs.append(graph)
        outs.append(res)
        pool = pool or graph.pool()
    for turn in range(3):
        for graph, (name, leaves, call), res in zip(graphs, calls, outs):
            out = call(*leaves)
            want = (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(res, want):
                assert torch.equal(x, y), (name, turn)


def test_bad_sizes_of_a_plan_raise():
    """What the C entries refuse by themselves comes back as an error, not as a launch."""
    from smsgate_amd import ops

    lib = ops.load_library()
    import ctypes

    plan = (ctypes.c_int * 6)()
    assert lib.sg_loss_plan(0, 5, 8, plan) and lib.sg_loss_plan(5, 5, 12, plan) and lib.sg_loss_plan(5, 0, 8, plan)
    assert lib.sg_attn_fwd(None, None, None, None, None, None, None, (ctypes.c_long * 9)(), 1, 5, 3, 2, 64, 1, 0, 1.0,
                           None) == 1
    assert lib.sg_embed_fwd(None, None, 1, None, None, 0, 5, 8, 1.0, 0, 1, None) == 1
