"""The training operators' autograd functions (ops/csrc/train_autograd.cpp): what autograd's
modes ask of them."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

dev = "cuda"


def _calls():
    from smsgate_amd.models import train_ops

    g = torch.Generator(device=dev).manual_seed(11)

    def normal(*s):
        return torch.randn(*s, generator=g, device=dev)

    ids = torch.randint(0, 500, (4, 60), generator=g, device=dev)
    add = torch.randint(-1, 500, (4, 60), generator=g, device=dev)
    labels = torch.randint(-1, 500, (4, 60), generator=g, device=dev)
    lengths = torch.tensor([60, 17], dtype=torch.int32, device=dev)
    return [
        ("embed", [normal(500, 64).requires_grad_()], lambda t: train_ops.embed_lookup(ids, t, add, scale=8.0)),
        ("attention", [normal(2, h, 60, 64).bfloat16().requires_grad_() for h in (4, 2, 2)],
         lambda q, k, v: train_ops.tiled_attention(q, k, v, lengths=lengths)),
        ("loss", [normal(4, 60, 64).half().requires_grad_(), normal(500, 64).half().requires_grad_()],
         lambda h, t: train_ops.lm_loss(h, t, labels, ignore_index=-1)),
    ]


def test_without_gradients_the_result_is_the_same():
    for name, leaves, call in _calls():
        a = call(*leaves)
        with torch.no_grad():
            b = call(*leaves)
        c = call(*(t.detach() for t in leaves))
        assert a.requires_grad and not b.requires_grad and not c.requires_grad, name
        assert torch.equal(a, b) and torch.equal(a, c), name


def test_each_input_alone():
    """Only one input asks for a gradient: the same bits as with all of them."""
    for name, leaves, call in _calls():
        out = call(*leaves)
        g = torch.ones_like(out)
        want = torch.autograd.grad(out, leaves, g)
        for i, w in enumerate(want):
            some = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
            (x,) = torch.autograd.grad(call(*some), some[i], g)
            assert torch.equal(x, w), (name, i)


def test_recomputed_in_the_backward():
    """Under checkpointing the forward runs again in autograd's thread, through its hooks."""
    for name, leaves, call in _calls():
        out = call(*leaves)
        g = torch.ones_like(out)
        want = torch.autograd.grad(out, leaves, g)
        again = checkpoint(call, *leaves, use_reentrant=False)
        assert torch.equal(out, again), name
        for x, w in zip(torch.autograd.grad(again, leaves, g), want):
            assert torch.equal(x, w), name


def test_in_place_changes_before_the_backward_are_seen():
    from smsgate_amd.models import train_ops

    q, k, v = (torch.randn(1, 2, 40, 64, device=dev).bfloat16() for _ in range(3))
    leaf = q.clone().requires_grad_()
    mid = leaf * 1
    out = train_ops.tiled_attention(mid, k, v)
    mid.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()


def test_a_penalty_on_gradients_raises():
    """Where a second derivative would be left out, there is an error instead."""
    for name, leaves, call in _calls():
        if name == "embed":
            continue  # linear: its gradient does not depend on the table
        out = call(*leaves).float().pow(2).sum()
        grads = torch.autograd.grad(out, leaves, create_graph=True)
        with pytest.raises(RuntimeError, match="again"):
            (out + sum(g.float().pow(2).sum() for g in grads)).backward()


def test_freed_after_the_backward():
    for name, leaves, call in _calls():
        out = call(*leaves)
        g = torch.ones_like(out)
        torch.autograd.grad(out, leaves, g)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(out, leaves, g)


def test_memory_goes_with_the_results():
    """Nothing outlives the call's tensors."""
    for name, leaves, call in _calls():
        for _ in range(2):
            out = call(*leaves)
            torch.autograd.grad(out, leaves, torch.ones_like(out))
            del out
            torch.cuda.synchronize()
            held = torch.cuda.memory_allocated()
            if _ == 0:
                first = held
        assert held == first, name


def test_capture_beside_a_living_eager_graph_is_refused():
    """The captured backward would end the process; the captured forward raises instead."""
    for name, leaves, call in _calls():
        alive = call(*leaves)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(graph):
                call(*leaves)
        want = torch.autograd.grad(alive, leaves, torch.ones_like(alive))
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*leaves)
            got = torch.autograd.grad(out, leaves, torch.ones_like(out))
            del out
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            for x, w in zip(got, want):
                assert torch.equal(x, w), name
