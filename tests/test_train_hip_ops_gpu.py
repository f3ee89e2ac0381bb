"""The training step with the embedding, attention and loss of this package
(TrainConfig.hip_ops): embed_lookup -> layers with tiled_attention -> lm_loss, as
train_extractor runs them together."""
import dataclasses

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

dev = "cuda"


def _rel(a, b):
    return float((a.float() - b.float()).norm() / (b.float().norm() + 1e-12))


def _weights(name="smollm-135m", layers=3, vocab=1024):
    from smsgate_amd.models.extractor import CONFIGS, ExtractorWeights

    cfg = dataclasses.replace(CONFIGS[name], layers=layers, vocab=vocab)
    return ExtractorWeights(cfg, device=dev, dtype=torch.float32, seed=5)


def _grads(w, loss):
    loss.backward()
    g = {n: p.grad.detach().clone() for n, p in w.named_parameters()}
    w.zero_grad(set_to_none=True)
    return g


@pytest.mark.parametrize("name", ["smollm-135m", "small", "smollm-360m"])
def test_step_matches_reference_forward(name):
    """Loss and every gradient of a padded batch against reference_forward with
    cross_entropy, both bf16 autocast over fp32 masters (the tolerances of
    tests/test_train_ops_gpu.py, whose forward this is)."""
    from smsgate_amd.models import train_ops
    from smsgate_amd.models.extractor import reference_forward

    w = _weights(name)
    g = torch.Generator(device=dev).manual_seed(3)
    B, T = 5, 77
    lens = torch.tensor([77, 40, 3, 64, 65], device=dev)
    ids = torch.randint(0, w.cfg.vocab, (B, T), generator=g, device=dev)
    add = torch.where(torch.rand(B, T, generator=g, device=dev) < 0.5,
                      torch.randint(0, w.cfg.vocab, (B, T), generator=g, device=dev), -1)
    labels = torch.randint(0, w.cfg.vocab, (B, T), generator=g, device=dev)
    labels[(torch.rand(B, T, generator=g, device=dev) < 0.6) | (torch.arange(T, device=dev) >= lens[:, None])] = -100
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        h = train_ops.fused_forward(w, ids, add, hip_ops=True, lengths=lens.int())
        loss = train_ops.lm_loss(h, w.embed.to(h.dtype), labels)
    got = _grads(w, loss)
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        hr = reference_forward(w, ids, compute_dtype=torch.float32, return_hidden=True, add_ids=add)
        sel = labels >= 0
        ref = F.cross_entropy((hr[sel] @ w.embed.t()).float(), labels[sel])
    want = _grads(w, ref)
    assert abs(float(loss) - float(ref)) <= 2e-2 * abs(float(ref))
    for b, n in enumerate(lens.tolist()):
        assert _rel(h[b, :n].detach(), hr[b, :n].detach()) < 2e-2
    for n in want:
        assert _rel(got[n], want[n]) < 5e-2, n


def test_lengths_change_no_labelled_row():
    """With and without lengths: the same bits in every row inside its sequence."""
    from smsgate_amd.models import train_ops

    w = _weights(layers=2)
    ids = torch.randint(0, w.cfg.vocab, (4, 70), device=dev)
    lens = torch.tensor([70, 33, 1, 64], dtype=torch.int32, device=dev)
    with torch.no_grad(), torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        a = train_ops.fused_forward(w, ids, hip_ops=True)
        b = train_ops.fused_forward(w, ids, hip_ops=True, lengths=lens)
        for i, n in enumerate(lens.tolist()):
            assert torch.equal(a[i, :n], b[i, :n])
        with pytest.raises(ValueError, match="hip_ops"):
            train_ops.fused_forward(w, ids, lengths=lens)


@pytest.mark.parametrize("fmt", ["qa", "span", "copy"])
def test_train_extractor_runs(fmt):
    """A few steps of each answer format through train_extractor: finite weights, and the
    same weights from the same seed (every sum of the new operators has a fixed order)."""
    from smsgate_amd.models.train import TrainConfig, train_extractor

    cfg = TrainConfig(model="small", steps=6, batch=16, n_examples=200, warmup=2, log_every=0, answer_format=fmt,
                      hip_ops=True, ema=0.0)
    a, b = (train_extractor(cfg, device="cuda", log=lambda *_: None) for _ in range(2))
    for (n, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert torch.isfinite(p).all(), n
        if fmt != "qa":  # the qa loss itself gathers by torch's atomics
            assert _rel(p, q) <= 1e-2, n
